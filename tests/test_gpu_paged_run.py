"""GPU: the paged operators as a program runs them: prompts packed and stored,
then steps of plan, store and tree attention in one captured graph, replayed
while the requests grow; every row against the plain implementation over the
request's own keys and values."""
import numpy as np
import pytest
import torch

from iris_amd import native, paged, scalars
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def dev(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


@pytest.mark.parametrize("heads, kv_heads, hd, window, scaled, page", [
    (8, 2, 64, 0, True, 16), (4, 1, 128, 40, False, 4), (6, 3, 80, 0, True, 32), (2, 1, 256, 70, False, 8)])
@pytest.mark.parametrize("captured", [False, True])
def test_prompts_then_steps(heads, kv_heads, hd, window, scaled, page, captured):
    rng = np.random.default_rng(hd + page)
    prompts, nodes, steps = [33, 1, 70, 16], 3, 6
    n, rows, kvw, qw = len(prompts), sum(prompts), kv_heads * hd, heads * hd
    parents = [-1, 0, 0]  # the token, and two drafts of what follows it: the second is kept
    scale = scalars.attention_scale_q32(hd) if scaled else 0
    stride = -(-(max(prompts) + 2 * steps + nodes) // page)
    pages = sum(-(-(p + 2 * steps + nodes) // page) for p in prompts) + 1
    draw = lambda *shape: (rng.normal(0, 65536, shape)).round().astype(np.int32)
    k_pages = torch.full((pages, kv_heads, page, hd), 99, dtype=torch.int32, device="cuda")
    v_pages = torch.full_like(k_pages, 98)
    cache = paged.PagedKv(k=k_pages.data_ptr(), v=v_pages.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    t = dict(lengths=dev([0] * n), added=dev(prompts), held=dev([0] * n), table=dev(np.full((n, stride), -1)),
             ring=dev(rng.permutation(pages)), ring_state=dev([0, pages]), row_start=dev([0] * (n + 1)), slots=dev([0] * rows),
             positions=dev([0] * rows), status=dev([0]))
    plan = paged.PagedPlan(**{x: y.data_ptr() for x, y in t.items()}, held_out=t["held"].data_ptr(),
                           ring_state_out=t["ring_state"].data_ptr(), requests=n, table_stride=stride, pages=pages,
                           page_size=page, max_rows=rows)
    q, k, v = draw(rows, qw), draw(rows, kvw), draw(rows, kvw)
    tq, tk, tv = dev(q), dev(k), dev(v)
    out = torch.zeros((rows, qw), dtype=torch.int32, device="cuda")
    packed = paged.PackedAttention(q=tq.data_ptr(), k=tk.data_ptr(), v=tv.data_ptr(), out=out.data_ptr(),
                                   row_start=t["row_start"].data_ptr(), q_stride=qw, k_stride=kvw, v_stride=kvw, out_stride=qw,
                                   sequences=n, rows=rows, max_length=max(prompts), heads=heads, kv_heads=kv_heads, head_dim=hd,
                                   window=window, scaled=int(scaled), scale_q32=scale)
    space = torch.empty(max(paged.packed_workspace_bytes(packed), 16), dtype=torch.uint8, device="cuda")
    paged.plan(plan)
    paged.store(cache, tk.data_ptr(), kvw, tv.data_ptr(), kvw, t["slots"].data_ptr(), rows)
    paged.attend_packed(packed, space.data_ptr(), space.numel())
    torch.cuda.synchronize()
    starts = np.concatenate([[0], np.cumsum(prompts)]).tolist()
    want = ref.packed(q, k, v, starts, heads, kv_heads, hd, window, scale, np.zeros((rows, qw), np.int32))
    assert t["status"].item() == 0 and np.array_equal(out.cpu().numpy(), want)
    keys = [k[a:b] for a, b in zip(starts[:-1], starts[1:])]
    vals = [v[a:b] for a, b in zip(starts[:-1], starts[1:])]

    # Steps: three rows a request.
    m = n * nodes
    sq, sk, sv = (torch.zeros((m, w), dtype=torch.int32, device="cuda") for w in (qw, kvw, kvw))
    step_out = torch.zeros((m, qw), dtype=torch.int32, device="cuda")
    t["parents"] = dev(parents * n)
    plan.parents, plan.max_rows = t["parents"].data_ptr(), m
    tree = paged.TreeAttention(q=sq.data_ptr(), out=step_out.data_ptr(), row_start=t["row_start"].data_ptr(),
                               lengths=t["lengths"].data_ptr(), parents=t["parents"].data_ptr(), table=t["table"].data_ptr(),
                               status=t["status"].data_ptr(), q_stride=qw, out_stride=qw, requests=n, rows=m, table_stride=stride,
                               max_nodes=nodes, max_positions=max(prompts) + 2 * steps + nodes, heads=heads, window=window,
                               scaled=int(scaled), scale_q32=scale)
    room = torch.empty(max(paged.tree_workspace_bytes(cache, tree), 16), dtype=torch.uint8, device="cuda")
    t["lengths"].copy_(dev(prompts))
    t["added"].fill_(nodes)
    # What is kept of a step, moved behind the last position by the next one's
    # store: the second draft's slot goes to the first's.
    kept_k, kept_v = torch.zeros_like(sk), torch.zeros_like(sv)

    def step(stream):
        paged.plan(plan, stream)
        paged.store(cache, sk.data_ptr(), kvw, sv.data_ptr(), kvw, t["slots"].data_ptr(), m, stream)
        paged.attend_tree(cache, tree, room.data_ptr(), room.numel(), stream)

    torch.cuda.synchronize()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(torch.cuda.current_stream().cuda_stream)
    for i in range(steps):
        q, k, v = draw(m, qw), draw(m, kvw), draw(m, kvw)
        for to, x in ((sq, q), (sk, k), (sv, v)):
            to.copy_(dev(x))
        if captured:
            g.replay()
        else:
            step(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert t["status"].item() == 0
        got, positions = step_out.cpu().numpy(), t["positions"].cpu().numpy()
        for b in range(n):
            length = len(keys[b])
            at = slice(b * nodes, b * nodes + nodes)
            assert positions[at].tolist() == [length, length + 1, length + 1]
            all_k, all_v = np.concatenate([keys[b], k[at]]), np.concatenate([vals[b], v[at]])
            seen, _ = ref.tree_mask(length, parents, window)
            for h in range(heads):
                c, kc = slice(h * hd, h * hd + hd), slice(h // (heads // kv_heads) * hd, (h // (heads // kv_heads) + 1) * hd)
                assert np.array_equal(got[at][:, c], ref.attend(q[at][:, c], all_k[:, kc], all_v[:, kc], seen, scale)), (i, b, h)
            # The token and its second draft are kept.
            keep = [b * nodes, b * nodes + 2]
            keys[b], vals[b] = np.concatenate([keys[b], k[keep]]), np.concatenate([vals[b], v[keep]])
        slots = t["slots"][:m].clone().view(n, nodes)
        kept_k.copy_(sk)
        kept_v.copy_(sv)
        slots[:, 0], slots[:, 2], slots[:, 1] = -1, slots[:, 1].clone(), -1
        moved = slots.reshape(-1).contiguous()
        paged.store(cache, kept_k.data_ptr(), kvw, kept_v.data_ptr(), kvw, moved.data_ptr(), m,
                    torch.cuda.current_stream().cuda_stream)
        t["lengths"] += 2
    torch.cuda.synchronize()
