"""GPU test of a decoder's step of several sequences as the documents have it: their code is what runs."""
import math
import os
import textwrap

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


def blocks():
    """The guide's two: the prompts and their indexes, a step.  And the step of the module's own text."""
    from cuvs_b200 import kv_cache
    with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
        text = f.read()
    text = text[text.index("**A decoder's step over a long context**"):]
    found = [part.split("```")[0] for part in text.split("```python\n")[1:3]]
    doc = kv_cache.__doc__
    doc = doc[doc.index("is::") + 4:doc.index("An index that several")]
    return found[0], found[1], "from cuvs_b200 import ivf_pq, kv_cache\nimport torch\n" + textwrap.dedent(doc)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k,n_probes", [(40, 4), (501, 8)])
def test_the_documented_step(dtype, k, n_probes):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cuvs_b200 import ivf_pq
    g = torch.Generator(device="cuda").manual_seed(7)
    prompts, n_heads, group, dim, window, page = [1500, 700, 2100], 2, 3, 64, 200, 64
    n_sequences, total = len(prompts), sum(prompts)

    def rows(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    width = max(prompts) // page + 1
    has = {"dtype": dtype, "n_pages": n_sequences * width, "n_heads": n_heads, "dim": dim, "n_sequences": n_sequences, "n_lists": 8,
           "window": window, "k": k, "params": ivf_pq.SearchParams(n_probes=n_probes),
           "pages": torch.randperm(n_sequences * width, generator=g, device="cuda").int().view(n_sequences, width),
           "prompt_keys": rows(total, n_heads, dim), "prompt_values": rows(total, n_heads, dim),
           "prompt_sequences": ints([i for i, n in enumerate(prompts) for _ in range(n)]),
           "prompt_positions": ints([p for n in prompts for p in range(n)]), "positions": ints(prompts), "lengths": ints([n + 1 for n in prompts]),
           "new_keys": rows(n_sequences, n_heads, dim), "new_values": rows(n_sequences, n_heads, dim),
           "queries": rows(n_sequences, n_heads * group, dim),
           "frequencies": torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64, device="cuda")}
    prompt, step, own_step = blocks()
    exec(prompt, has)
    exec(own_step, has)
    before = has["out"].clone(), has["lse"].clone(), has["candidates"].clone()
    exec(step, has)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (has["out"], has["lse"], has["candidates"])))

    keys, values, q = (has[name].double() for name in ("keys", "values", "q"))
    pages, scale = has["pages"].long(), dim ** -0.5
    for i, n in enumerate(prompts):
        at = torch.arange(n + 1, device="cuda")
        own_slots = pages[i, at // page] * page + at % page
        for j in range(n_heads * group):
            named = has["candidates"][i, j]
            named = named[(named >= 0) & (named < n_sequences * width * page)]
            far = own_slots[:n + 1 - window]
            assert torch.isin(named, far).all() and named.unique().numel() == named.numel()     # its own, and none of the window
            assert named.numel() == min(k, far.numel()) or n_probes < 8
            slots = torch.cat((own_slots[n + 1 - window:], named))
            key, value = (t[slots // page, slots % page, j // group] for t in (keys, values))
            scores = scale * (key @ q[i, j])
            lse = torch.logsumexp(scores, 0)
            p = torch.exp(scores - lse)
            # as two 32-bit softmaxes, whose parts are rounded to their type and then joined and rounded once more
            total = 2 * (dim + 4) * U * scale * (key.abs() @ q[i, j].abs()).max() + 2.0 ** -20 + (slots.numel() + 600) * U
            parts = torch.stack((has["near"][i, j], has["far"][i, j])).double().abs().amax(0)
            tol = 2 * total * (p @ value.abs()).max() + torch.finfo(dtype).eps / 2 * (parts + (p @ value).abs()) + 2.0 ** -24
            assert ((has["out"][i, j].double() - p @ value).abs() <= tol).all(), (i, j)
            assert abs(has["lse"][i, j].item() - lse.item()) <= total + 4 * U * (1 + abs(lse.item()))
            if named.numel() == far.numel():
                assert math.isclose(lse.item(), torch.logsumexp(scale * (keys[own_slots // page, own_slots % page, j // group] @ q[i, j]), 0).item(),
                                    rel_tol=1e-9)                                               # every far key was found: attention to all
