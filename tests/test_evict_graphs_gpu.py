"""Trees, sums of weights, selection and moving of tokens captured into graphs, replayed with new inputs, on streams of their own, and in
pools of more than 2^32 bytes: the same answers as plain calls (the kernels have a fixed order of operations, so bit for bit)."""
import pytest
import torch

from leankv_b200 import attention, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, H, GRP, D, P, PER = 2, 2, 4, 128, 16, 40


def _inputs(seed, n, kind=8):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(lens=torch.tensor([600, 411], dtype=torch.int32, device=DEV))
    s["table"] = torch.randperm(B * PER, generator=torch.Generator().manual_seed(seed)).view(B, PER).to(torch.int32).to(DEV)
    for t in "kv":
        if kind == 8:
            s[t] = torch.randint(-127, 128, (B * PER, H, P, D), dtype=torch.int8, device=DEV, generator=g)
            s[t + "s"] = torch.exp(torch.randn(B * PER, H, P // 16, device=DEV, generator=g)) / 100
        else:
            s[t] = ops.quantize(torch.randn(B * PER, H, P, D, device=DEV, generator=g), kind if t == "k" else 4)
            s[t + "s"] = None
    s["q"] = torch.randn(B, H * GRP, n, D, device=DEV, generator=g).bfloat16()
    s["lse"] = 5 + torch.rand(B, H * GRP, n, device=DEV, generator=g)
    s["w"] = torch.rand(B * PER, H, P, device=DEV, generator=g)
    i = torch.arange(n, device=DEV)
    s["parents"] = ((torch.rand(B, n, device=DEV, generator=g) * (i + 1)).long() - 1).to(torch.int32)
    return s


def _tree(s):
    return attention.attention_q8_paged(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"], tree=ops.draft_tree(s["parents"]))


def _weights(s):
    return attention.attention_weights_paged(s["q"], s["k"], s["table"], s["lens"], s["lse"], s["w"], k_scale=s["ks"], decay=0.5)


def _select(s):
    return ops.select_tokens(s["w"], s["table"], s["lens"], 300, sinks=4, recent=16)


def _evict(s):
    ops.kv_move_paged(s["k"], s["v"], s["table"], _select(s), k_scale=s["ks"], v_scale=s["vs"], weights=s["w"])
    return [s[t] for t in ("k", "v", "ks", "vs", "w") if s[t] is not None]


CALLS = [(_tree, 5, 8), (_tree, 30, 8), (_tree, 150, 8), (_weights, 1, 8), (_weights, 6, 8), (_weights, 90, 8), (_weights, 1, 3), (_select, 1, 8),
         (_evict, 1, 8), (_evict, 1, 3)]


def _list(x):
    return [t.clone() for t in (x if isinstance(x, list) else [x])]


@pytest.mark.parametrize("call,n,kind", CALLS)
def test_captured_and_replayed_with_new_inputs(call, n, kind):
    state = _inputs(1, n, kind)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(_inputs(2, n, kind))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(state)
    for seed in (3, 4):
        fresh = _inputs(seed, n, kind)
        want = _list(call(_inputs(seed, n, kind)))
        for k, t in state.items():
            if t is not None:
                t.copy_(fresh[k])
        graph.replay()
        for a, b in zip(_list(out), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("call,n,kind", CALLS)
def test_calls_that_overlap_on_two_streams(call, n, kind):
    states = [_inputs(s, n, kind) for s in (5, 6)]
    want = [_list(call(_inputs(s, n, kind))) for s in (5, 6)]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    got = []
    for state, stream in zip(states, streams):
        with torch.cuda.stream(stream):
            got.append(call(state))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(_list(g), w):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", [8, 4])
def test_pools_of_more_than_2_to_the_32_bytes(kind):
    """Pages at the end of pools of 2^32 bytes and more."""
    page_bytes = H * P * (D if kind == 8 else 72)
    pages = (1 << 32) // page_bytes + 200
    small, far = _inputs(7, 40 if kind == 8 else 1, kind), _inputs(7, 40 if kind == 8 else 1, kind)
    for t in ("k", "v", "ks", "vs", "w"):
        if far[t] is not None:
            big = torch.zeros(pages, *far[t].shape[1:], dtype=far[t].dtype, device=DEV)
            big[-B * PER:] = far[t]
            far[t] = big
    far["table"] = far["table"] + (pages - B * PER)
    for call in ([_tree] if kind == 8 else []) + [_weights, _select, _evict]:
        a, b = call(small), call(far)
        for x, y in zip(_list(a), [t[-B * PER:] if t.shape[0] == pages else t for t in (b if isinstance(b, list) else [b])]):
            assert torch.equal(x, y)
