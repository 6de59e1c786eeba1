"""Beam search over a 4-bit KV cache that is kept to a token budget.

A toy attention model (random weights) generates with every cache operator in the order a
serving loop calls them:

  prompt   kv4_append of the prompt's K and V, one fork per beam (blocks shared)
  step     kv4_append of each beam's new token, kv4_paged_attn_decode with accumulated
           weights, beam_select over the logits, beam_gather of the token histories, weights
           and positions, reorder_sequences of the block tables
  budget   when a beam's cache passes budget + slack: cow_blocks (its blocks become its own),
           evict_tokens per layer, truncate_sequence

Run:  python examples/evicting_beams.py [--steps 96] [--beams 4] [--budget 96]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from lattice_b200 import CacheFormat, kcmm, make_config  # noqa: E402
from lattice_b200.workloads import library  # noqa: E402

LAYERS, HQ, HKV, D, VOCAB, BS = 2, 8, 2, 64, 1000, 16


class Toy:
    """x -> x + attention(x) per layer, tied embedding; positions enter through K alone."""

    def __init__(self, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        hidden = HQ * D
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.embed = r(VOCAB, hidden) * 0.5
        self.wq, self.wk, self.wv = ([r(hidden, n) * hidden ** -0.5 for _ in range(LAYERS)]
                                     for n in (HQ * D, HKV * D, HKV * D))
        self.pos = r(1 << 14, HKV * D) * 0.3

    def kv(self, layer, x, position):
        k = x @ self.wk[layer] + self.pos[position]
        return k.bfloat16().contiguous(), (x @ self.wv[layer]).bfloat16().contiguous()


def generate(steps: int = 96, beams: int = 4, prompt: int = 70, budget: int = 96, sinks: int = 4,
             recent: int = 32, slack: int = 16, seed: int = 0) -> dict:
    torch.cuda.set_device(0)
    model, stream = Toy(seed), torch.cuda.current_stream().cuda_stream
    # a beam holds at most max(prompt, budget + slack) + 1 tokens at a time
    most = max(prompt, budget + slack) + BS
    pool = library().create_pool(make_config(
        num_layers=LAYERS, kv_heads=HKV, head_dim=kcmm.kv4_row_elems(D), max_batch=3 * beams,
        max_seq_len=-(-most // BS) * BS, block_size=BS))
    tables = kcmm.StepTables(pool, beams)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    try:
        def append(layer, seqs, positions, x, position):
            """K and V of one token a sequence (or of the whole prompt) into their slots."""
            slots = [pool.block_table(s)[p // BS] * BS + p % BS for s, p in zip(seqs, positions)]
            d_slots = torch.tensor(slots, device="cuda")
            k, v = model.kv(layer, x, position)
            pool.kv4_append(layer, slot_mapping_ptr=d_slots.data_ptr(),
                            block_offsets_f16_ptr=tables.block_offsets_ptr,
                            block_offsets_f16_len=pool.total_blocks(), num_tokens=len(slots),
                            head_dim=D, k_src_ptr=k.data_ptr(), v_src_ptr=v.data_ptr(),
                            stream_ptr=stream)

        def grow(seq, tokens):
            while len(pool.block_table(seq)) * BS < tokens:
                pool.append_block_to_sequence(seq, pool.alloc_blocks(1)[0])
            pool.update_seq_len(seq, tokens)

        # prompt: cached once, then shared by the beams
        first = pool.register_sequence(pool.alloc_blocks(-(-prompt // BS)))
        pool.update_seq_len(first, prompt)
        tables.sync([first], stream)
        ids = torch.arange(prompt, device="cuda") * 7 % VOCAB
        for layer in range(LAYERS):
            append(layer, [first] * prompt, range(prompt), model.embed[ids],
                   torch.arange(prompt, device="cuda"))
        seqs = [first] + [pool.fork_sequence(first) for _ in range(beams - 1)]

        stride, length, position = most, prompt, prompt
        weights = [torch.zeros(2, beams, HKV, stride, device="cuda") for _ in range(LAYERS)]
        places = [i32(2, beams, HKV, stride) for _ in range(LAYERS)]  # stored positions
        history, kept = i32(2, beams, steps), i32(beams)
        scores = torch.full((1, beams), -float("inf"), device="cuda")
        scores[0, 0] = 0.0  # the beams start equal: only the first counts
        new_scores, parents, tokens = torch.empty_like(scores), i32(1, beams), i32(1, beams)
        new_lens, token = i32(beams), ids[-1].repeat(beams)
        cur, cuts = 0, 0
        # the prompt's last blocks are written next: beams that share them get their own
        for step in range(steps):
            shared = [(s, length // BS) for s in seqs
                      if length // BS < len(pool.block_table(s))
                      and pool.refcount(pool.block_table(s)[length // BS]) > 1]
            if shared:
                pool.cow_blocks([s for s, _ in shared], [b for _, b in shared], stream)
            for s in seqs:
                grow(s, length + 1)
            tables.sync(seqs, stream)
            x = model.embed[token.long()]
            for layer in range(LAYERS):
                append(layer, seqs, [length] * beams, x,
                       torch.full((beams,), position, device="cuda"))
                q = (x @ model.wq[layer]).bfloat16().view(beams, HQ, D).contiguous()
                out, w = torch.empty_like(q), weights[layer][cur]
                pool.kv4_paged_attn_decode(
                    layer, query_ptr=q.data_ptr(), out_ptr=out.data_ptr(),
                    block_tables_ptr=tables.block_tables_ptr, seq_lens_ptr=tables.seq_lens_ptr,
                    block_offsets_f16_ptr=tables.block_offsets_ptr, batch=beams, num_q_heads=HQ,
                    kv_heads=HKV, head_dim=D, block_size=BS,
                    max_blocks_per_seq=-(-most // BS), scale=D ** -0.5,
                    weights_in_ptr=w.data_ptr(), weights_out_ptr=w.data_ptr(),
                    weights_row_stride=stride, stream_ptr=stream)
                x = x + out.float().view(beams, -1)
            length, position = length + 1, position + 1

            logits = (x @ model.embed.T * 0.02).contiguous()
            pool.beam_select(logits_ptr=logits.data_ptr(), dtype="f32",
                             scores_in_ptr=scores.data_ptr(), batch=1, beams=beams, vocab=VOCAB,
                             n_select=beams, scores_out_ptr=new_scores.data_ptr(),
                             parents_out_ptr=parents.data_ptr(),
                             tokens_out_ptr=tokens.data_ptr(), stream_ptr=stream)

            def gather(buf, **kw):
                pool.beam_gather(src_ptr=buf[cur].data_ptr(), dst_ptr=buf[1 - cur].data_ptr(),
                                 row_bytes=buf[0, 0].numel() * 4, parents_ptr=parents.data_ptr(),
                                 batch=1, beams=beams, n_select=beams, stream_ptr=stream, **kw)
            gather(history, tokens_ptr=tokens.data_ptr(), token_index=step)
            for layer in range(LAYERS):
                gather(weights[layer])
                gather(places[layer])
            cur = 1 - cur
            pool.reorder_sequences(seqs, parents[0].tolist(), stream)
            scores, new_scores = new_scores, scores
            token = tokens[0].clone()

            if length > budget + slack:
                pairs = [(s, b) for s in seqs for b in range(-(-budget // BS))]
                pool.cow_blocks([s for s, _ in pairs], [b for _, b in pairs], stream)
                tables.sync(seqs, stream)
                nxt = torch.full((beams,), position, dtype=torch.int32, device="cuda")
                for layer in range(LAYERS):
                    w, p = weights[layer][cur], places[layer][cur]
                    pool.evict_tokens(
                        layer, cache_format=CacheFormat.KV4, head_dim=D,
                        block_tables_ptr=tables.block_tables_ptr,
                        seq_lens_ptr=tables.seq_lens_ptr,
                        block_offsets_f16_ptr=tables.block_offsets_ptr, batch=beams,
                        max_blocks_per_seq=-(-most // BS), budget=budget, sinks=sinks,
                        recent=recent, weights_in_ptr=w.data_ptr(), weights_out_ptr=w.data_ptr(),
                        weights_row_stride=stride, positions_in_ptr=p.data_ptr(),
                        positions_out_ptr=p.data_ptr(), next_positions_ptr=nxt.data_ptr(),
                        kept_lens_ptr=kept.data_ptr(), new_lens_ptr=new_lens.data_ptr(),
                        stream_ptr=stream)
                for s in seqs:
                    pool.truncate_sequence(s, budget)
                kept.fill_(budget)
                length, cuts = budget, cuts + 1
        torch.cuda.synchronize()
        status = pool.kernel_status()
        return {"tokens": history[cur].cpu(), "scores": scores[0].cpu(), "cuts": cuts,
                "cached": length, "positions": places[0][cur][:, :, :int(kept[0])].cpu(),
                "position": position, "blocks": pool.blocks_in_use(), "kernel_status": status,
                "block_tables": [pool.block_table(s) for s in seqs]}
    finally:
        tables.destroy()
        pool.destroy()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=96)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--budget", type=int, default=96)
    a = ap.parse_args()
    r = generate(steps=a.steps, beams=a.beams, budget=a.budget)
    for s, t in zip(r["scores"].tolist(), r["tokens"].tolist()):
        print(f"{s:9.3f}  {' '.join(map(str, t[:12]))} ...")
    print(f"{r['position']} positions seen, {r['cached']} cached after {r['cuts']} evictions, "
          f"{r['blocks']} blocks in use")


if __name__ == "__main__":
    main()
