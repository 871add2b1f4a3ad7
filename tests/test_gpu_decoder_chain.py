"""A decode loop that stays on the device: prompts, then steps replayed from one CUDA graph. Each step takes the
embedding rows of the last drawn ids through two attention layers (cuBLAS products standing in for the rest of
the model, ssb_norm_rope_append and ssb_attend_rows for their middle) to logits, draws the next ids and
gathers their rows (ssb_sample_embed_rows); the lengths grow on the device and nothing is read back between
steps. After every step each layer's new cache slots, query rows and attention rows are checked against the
plain forms in 64 bits on what the layer was given, the draws against the logits, and the fused LM head against
the draws."""
import pytest

import decoder_plain as plain
import speech_sampler as ss

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, VOCAB, PAGE = 8, 4, 64, 512, 2048, 16


def layer_weights(torch, g):
    width = (HEADS + 2 * KV) * DIM
    return dict(qkv=(torch.randn(HIDDEN, width, device="cuda", generator=g) / HIDDEN ** 0.5).to(torch.bfloat16),
                out=(torch.randn(HEADS * DIM, HIDDEN, device="cuda", generator=g) / HIDDEN ** 0.5).to(torch.bfloat16),
                q_weight=1 + 0.2 * torch.randn(DIM, device="cuda", generator=g),
                k_weight=1 + 0.2 * torch.randn(DIM, device="cuda", generator=g))


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_prompts_then_captured_steps(engine, window, sinks):
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    prompts, steps = [37, 1, 130], 7
    lens = [n + steps for n in prompts]
    layers = [layer_weights(torch, g) for _ in range(2)]
    cases = [plain.Case(lens, [1, 1, 1], HEADS, KV, DIM, torch.bfloat16, PAGE, seed=i, fill=float("nan")) for i in range(2)]
    for c in cases:
        c.table = cases[0].table  # one page table for all layers
        c.k.fill_(float("nan")), c.v.fill_(float("nan"))  # nothing is there yet
    caches = [c.cache() for c in cases]
    embedding = torch.randn(VOCAB, HIDDEN, device="cuda", generator=g).to(torch.bfloat16)
    inv_freq = 1e4 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") / (DIM // 2))
    length = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    scale = DIM ** -0.5

    def run_layers(x, record, **rows):
        n = x.shape[0]
        for i, w in enumerate(layers):
            qkv = x @ w["qkv"]
            q, k, v = (p.view(n, -1, DIM) for p in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
            stream = torch.cuda.current_stream()
            q_out = engine.norm_rope_append(q, k, v, caches[i], length, inv_freq, w["q_weight"], w["k_weight"], 1e-6,
                                            q_out=record[i]["q"], stream=stream, **rows)
            engine.attend(q_out, caches[i], length, scale, window, sinks, max_length=max(lens), out=record[i]["out"],
                          stream=stream, **rows)
            record[i]["qkv"].copy_(qkv)
            x = x + record[i]["out"].flatten(1) @ w["out"]
        return x

    def buffers(n):
        return [dict(q=torch.empty(n, HEADS, DIM, dtype=torch.bfloat16, device="cuda"),
                     out=torch.empty(n, HEADS, DIM, dtype=torch.bfloat16, device="cuda"),
                     qkv=torch.empty(n, (HEADS + 2 * KV) * DIM, dtype=torch.bfloat16, device="cuda")) for _ in layers]

    def check(record, rows, at):
        """Each layer's rows of this call: sequence s has rows[s] of them, up to position at[s]."""
        where = [(s, p) for s in range(3) for p in range(at[s] - rows[s], at[s])]
        positions = torch.tensor([p for _, p in where], device="cuda")
        page = torch.tensor([int(cases[0].table[s, p // PAGE]) for s, p in where], device="cuda")
        for c, w, r in zip(cases, layers, record):
            q, k, v = (p.view(len(where), -1, DIM) for p in r["qkv"].split([HEADS * DIM, KV * DIM, KV * DIM], 1))
            for x, weight, got in ((q, w["q_weight"], r["q"]), (k, w["k_weight"], c.k[page, positions % PAGE])):
                want, err = plain.norm_rope(x, weight, 1e-6, positions, inv_freq, False)
                assert torch.all((got.double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err))
            assert torch.equal(c.v[page, positions % PAGE], v)
            c.lens, c.rows, c.total, c.q = at, rows, len(where), r["q"]
            plain.check_attend(c, r["out"], None, scale, window, sinks)

    ids = torch.randint(0, VOCAB, (sum(prompts),), device="cuda", generator=g)
    row_start = torch.tensor([0, 37, 38, 168], dtype=torch.int32, device="cuda")
    record = buffers(sum(prompts))
    x = run_layers(embedding[ids], record, row_start=row_start, max_rows=max(prompts))
    torch.cuda.synchronize()
    check(record, prompts, prompts)

    hidden = x[row_start[1:].long() - 1].contiguous()
    logits = torch.empty(3, VOCAB, device="cuda")
    drawn, status = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    rows = torch.empty(3, HIDDEN, dtype=torch.bfloat16, device="cuda")
    fused = torch.empty(3, dtype=torch.int32, device="cuda")
    record = buffers(3)
    greedy = ss.params(greedy=True)

    def draw():
        torch.matmul(hidden.float(), embedding.float().T, out=logits)
        engine.sample_embed(logits, greedy, embedding, rows, ids=drawn, status=status, stream=torch.cuda.current_stream())
        engine.lm_head_argmax(hidden, embedding, fused, stream=torch.cuda.current_stream())

    def step():
        length.add_(1)
        hidden.copy_(run_layers(rows, record))
        draw()

    draw()
    kept = (rows.clone(), hidden.clone(), length.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # eager once, as graphs ask for
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for buffer, value in zip((rows, hidden, length), kept):
        buffer.copy_(value)
    for i in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        check(record, [1, 1, 1], [n + i + 1 for n in prompts])
        assert length.tolist() == [n + i + 1 for n in prompts] and status.tolist() == [ss.ROW_OK] * 3
        assert torch.equal(drawn.long(), logits.argmax(1)) and torch.equal(rows, embedding[drawn.long()])
        best = logits.topk(2, dim=1).values
        for r in range(3):  # the fused head sums in another order: within 1e-3 of a tie either may win
            assert int(fused[r]) == int(drawn[r]) or float(best[r, 0] - logits[r, int(fused[r])]) <= 1e-3
