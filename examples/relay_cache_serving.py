"""A serving loop on the 4-bit relay cache: a shared prompt, conversations that fork, grow and end.

    python examples/relay_cache_serving.py [--sequences 64] [--prefix 4096] [--steps 64]

One relay-attention layer of 16 heads of width 128.  The shared prompt is a row of the page table of its own, so
that its pages follow when the pool is compacted.  Every step reserves the next token's page (copying a page that
another conversation still shares), appends the token's key and value, and attends over [prompt ; own tokens].
At the end the last step is repeated by ``relay_merge_decode`` on the cache's values read back as dense tensors.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import delta_block_lm_b200 as dbl  # noqa: E402

H, D, PAGE = 16, 128, 64


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--sequences", type=int, default=64)
    ap.add_argument("--prefix", type=int, default=4096)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args(argv)
    dev, n = torch.device("cuda:0"), a.sequences
    torch.manual_seed(0)

    def tokens(*shape):  # keys and values of new tokens
        return [torch.randn(*shape, H, D, device=dev).to(torch.bfloat16) for _ in "kv"]

    ints = lambda x: torch.tensor(x, device=dev, dtype=torch.int32)  # noqa: E731
    longest = a.prompt + a.steps
    width = max(-(-longest // PAGE), -(-a.prefix // PAGE))
    pool = dbl.relay_cache_pool(n * (-(-longest // PAGE) + 1) + -(-a.prefix // PAGE), H, D, PAGE, device=dev)
    table = torch.full((n + 1, width), -1, device=dev, dtype=torch.int32)  # the last row: the shared prompt
    lengths = torch.zeros(n + 1, device=dev, dtype=torch.int32)
    refs = torch.zeros(len(pool), device=dev, dtype=torch.int32)

    def write(counts, k, v):
        nonlocal table, lengths, refs
        counts = ints(counts)
        table, refs, missing = dbl.relay_cache_reserve(pool, table, lengths, refs, counts)
        lengths = dbl.relay_cache_append(pool, table, lengths, k, v, counts=counts)
        return missing

    def attend(q):
        return dbl.relay_cache_attention(q, pool, table[:n], lengths[:n], prefix_pages=table[n], prefix_len=a.prefix)

    # the shared prompt, and the first half of the conversations
    half = max(1, n // 2)
    missing = write([0] * n + [a.prefix], *tokens(n + 1, a.prefix))
    missing = missing + write([a.prompt] * half + [0] * (n + 1 - half), *tokens(n + 1, a.prompt))
    # the other half continues from them and shares their pages until it writes
    table, lengths, refs = dbl.relay_cache_fork(pool, table, lengths, refs, ints(list(range(n - half))),
                                                ints(list(range(half, n))))
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(a.steps):
        if step == a.steps // 2:  # one conversation ends, another begins in its place; holes close
            table, lengths, refs = dbl.relay_cache_release(pool, table, lengths, refs, ints([0]))
            table, refs, used = dbl.relay_cache_compact(pool, table, refs)
        if step == 3:
            begin.record()
        missing = missing + write([1] * n + [0], *tokens(n + 1, 1))
        q = torch.randn(n, H, D, device=dev).to(torch.bfloat16)
        out, row_max, row_sum = attend(q)
    end.record()
    torch.cuda.synchronize()
    if missing.item():
        raise SystemExit(f"the pool lacked {missing.item()} pages")

    # the same attention on dense tensors
    own = int(lengths[:n].max())
    k, v = dbl.relay_cache_read(pool, table, lengths, tokens=max(own, a.prefix))
    dense = lambda x: x[:n, :own].transpose(1, 2).contiguous()  # noqa: E731
    shared = lambda x: x[n, :a.prefix].transpose(0, 1).contiguous()  # noqa: E731
    want, _, _ = dbl.relay_merge_decode(q, shared(k), shared(v), dense(k), dense(v), own_len=lengths[:n])
    err = float((out.float() - want.float()).norm() / want.float().norm())
    tokens_held = int(lengths.sum())
    print(f"{n} sequences, prompt {a.prefix} + {a.prompt}, {a.steps} steps: "
          f"{begin.elapsed_time(end) / max(1, a.steps - 3) * 1e3:.0f} us a step with its inputs")
    print(f"{tokens_held} tokens held, {int((refs > 0).sum())} pages in use ({int(used)} after compaction), "
          f"{int((refs > 0).sum()) * pool[0].numel() / 2 ** 20:.0f} MiB; dense bf16: "
          f"{tokens_held * H * D * 4 / 2 ** 20:.0f} MiB")
    print(f"relative difference to relay_merge_decode on the values read back: {err:.2e}")
    return err


if __name__ == "__main__":
    main()
