"""A long context in an 8-bit cache, cut down by attention weight: one attention layer's calls as a serving loop makes them.

A prompt goes into the cache in chunks (append + prefill). The last tokens' attention weights start a running sum per key
and kv head. Then rounds of drafts: append the drafts (they stay in the fp16 tail), attend, keep the accepted ones, add
the round's weights. When the cache holds more than the limit, the heaviest keys move into a smaller cache (the first and
the last tokens always stay) and the rounds go on there; new keys keep the RoPE rotation of their true position.

    python examples/long_context.py [--prompt 8192] [--rounds 40] [--limit 4096] [--budget 2048] [--format int8|e4m3]

Random K, V and queries stand in for a model's projections. Prints the memory and the time per round; needs a B200."""
import argparse
import pathlib
import sys

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "lfm3-1.7b-mi50_b200"))

import torch  # noqa: E402

import lfm3attn as la  # noqa: E402

Q_HEADS, KV_HEADS, HEAD_DIM, DRAFTS = 32, 8, 64, 8
SINK, RECENT = 4, 128


def run(prompt=8192, rounds=40, limit=4096, budget=2048, fmt="int8", chunk=2048, seed=0):
    """Returns what the loop did: tokens generated, evictions, the last output and the final cache."""
    mode = la.MODE_I8BLK if fmt == "int8" else la.MODE_E4M3BLK
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rows(n, heads):
        return torch.randn(n, heads, HEAD_DIM, generator=gen, device="cuda").half()

    positions = prompt + rounds * DRAFTS + DRAFTS
    rope = torch.from_numpy(la.rope_table(1e6, 1.0, HEAD_DIM, positions)).view(torch.float16).cuda()
    cache = la.LayerCache8(mode, KV_HEADS, HEAD_DIM, prompt + 128)
    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        cache.append(rows(n, KV_HEADS), rows(n, KV_HEADS), rope=rope)
        cache.prefill(rows(n, Q_HEADS), at)

    # The weights of the prompt's last tokens, and room for keys to come.
    m = min(32, prompt)
    q = rows(m, Q_HEADS)
    lse = torch.empty(m, Q_HEADS, device="cuda")
    cache.verify(q, cache.length - m, lse=lse)
    weights = torch.zeros(KV_HEADS, positions, device="cuda")
    cache.key_weights(q, lse, cache.length - m, out=weights)

    workspace = cache.workspace(DRAFTS, Q_HEADS)
    lse = torch.empty(DRAFTS, Q_HEADS, device="cuda")
    position, evictions, out = prompt, 0, None
    accepted = torch.randint(1, DRAFTS + 1, (rounds,), generator=torch.Generator().manual_seed(seed)).tolist()
    for keep_drafts in accepted:
        if cache.length > limit:
            smaller = la.LayerCache8(mode, KV_HEADS, HEAD_DIM, limit + 128)
            _, kept = cache.evict(weights, budget, SINK, RECENT, smaller)
            weights = torch.zeros(KV_HEADS, positions, device="cuda")
            weights[:, :budget] = kept
            cache, evictions = smaller, evictions + 1
            workspace = cache.workspace(DRAFTS, Q_HEADS)
        slot = cache.length
        # The cache's slots have moved on from the positions: the RoPE rows are those of the true positions.
        cache.append(rows(DRAFTS, KV_HEADS), rows(DRAFTS, KV_HEADS), rope=rope[position - slot:], draft=True)
        q = rows(DRAFTS, Q_HEADS)
        out = cache.verify(q, slot, lse=lse, workspace=workspace)
        cache.truncate(slot + keep_drafts)
        position += keep_drafts
        # The accepted tokens' weights on top of the sum so far (a little of it forgotten each round).
        cache.key_weights(q[:keep_drafts], lse[:keep_drafts], slot, prev=weights, decay=0.99, out=weights)
    la.sync()
    return {"position": position, "evictions": evictions, "out": out, "cache": cache, "weights": weights}


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--prompt", type=int, default=8192)
    p.add_argument("--rounds", type=int, default=40)
    p.add_argument("--limit", type=int, default=4096)
    p.add_argument("--budget", type=int, default=2048)
    p.add_argument("--format", choices=["int8", "e4m3"], default="int8")
    a = p.parse_args()
    if not SINK + RECENT <= a.budget <= a.limit:
        p.error("need %d <= budget <= limit" % (SINK + RECENT))
    run(a.prompt, 2, a.limit, a.budget, a.format)
    start, end = torch.cuda.Event(True), torch.cuda.Event(True)
    start.record()
    got = run(a.prompt, a.rounds, a.limit, a.budget, a.format)
    end.record()
    torch.cuda.synchronize()
    cache = got["cache"]
    print("%d tokens, %d evictions, %d in the cache (%.1f MB), %.2f ms in all" % (
        got["position"], got["evictions"], cache.length, (cache.pool.numel() + cache.tail.numel()) / 1e6,
        start.elapsed_time(end)))


if __name__ == "__main__":
    main()
