"""A paged cache of keys and values in plain torch (64 bits), for the tests of gptb200_kv_pages_* and gptb200_attention_paged."""
import torch

LOW, HIGH = -117, 119   # range of a row's power of two


def codes_of(x):
    """x [..., dim] in float64 -> (e4m3 codes' values in float64, exponents + 127 as uint8), from the definition: the smallest power of two whose 448-fold reaches the
    largest finite value, codes rounded to nearest even, what is not finite a NaN."""
    finite = torch.isfinite(x)
    y = torch.where(finite, x, torch.zeros_like(x))
    most = y.abs().amax(-1)
    e = torch.full_like(most, LOW).to(torch.int64)
    powers = torch.ldexp(torch.ones(HIGH - LOW + 1, dtype=torch.float64), torch.arange(LOW, HIGH + 1)).to(x.device)
    e = torch.searchsorted(448.0 * powers, most.contiguous()).clamp(max=HIGH - LOW) + LOW
    z = y / powers[e - LOW][..., None]
    size = torch.frexp(z.abs().clamp(min=2.0 ** -6))[1] - 1                 # exponent of the value, subnormals share the smallest normal's
    step = torch.ldexp(torch.ones_like(z), size - 3)
    code = (torch.round(z / step) * step).clamp(-448.0, 448.0)
    return torch.where(finite, code, torch.full_like(code, float("nan"))), (e + 127).to(torch.uint8)


class Cache:
    """Pages filled with other numbers (NaN where `poison`), tables of shuffled pages, and the three arrays of a call."""

    KINDS = {"bf16": 0, "f32": 1, "e4m3": 2}
    TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}

    def __init__(self, kind, lengths, counts, kv_heads, dim, page, seed=0, extra_rows=0, poison=False, spread=0.7, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.lengths, self.counts, self.kv_heads, self.dim, self.page = kind, list(lengths), list(counts), kv_heads, dim, page
        held = [-(-max(n, 0) // page) for n in lengths]
        self.num_pages = sum(held) + spare
        self.pitch = max(held + [0]) + 1
        order = torch.randperm(self.num_pages, generator=g).tolist()
        self.used = order[:sum(held)]
        table = torch.full((len(lengths), self.pitch), -1, dtype=torch.int32)   # what no row needs is no page's number
        at = 0
        for s, n in enumerate(held):
            table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table_cpu = table
        starts = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        starts[1:] = torch.tensor(self.counts, dtype=torch.int32).cumsum(0)
        self.starts_cpu, self.rows = starts, int(starts[-1]) + extra_rows
        x = torch.randn(self.num_pages, 2, kv_heads, page, dim, generator=g, dtype=torch.float64)
        x *= torch.exp(spread * torch.randn(self.num_pages, 2, kv_heads, page, 1, generator=g, dtype=torch.float64))
        if kind == "e4m3":
            codes, self.scales_cpu = codes_of(x)
            self.values = torch.ldexp(codes, self.scales_cpu[..., None].int() - 127)
            self.data_cpu = codes.to(torch.float32).to(torch.float8_e4m3fn)
        else:
            self.scales_cpu = None
            self.data_cpu = x.to(self.TYPES[kind])
            self.values = self.data_cpu.double()
        if poison:   # everything behind a sequence's last token, and pages that nobody has
            bad = torch.ones(self.num_pages, page, dtype=torch.bool)
            for s, n in enumerate(self.lengths):
                for i in range(max(n, 0)):
                    bad[int(table[s, i // page]), i % page] = False
            mask = bad[:, None, None, :, None].expand_as(self.values)
            self.data_cpu = self.data_cpu.float().masked_fill(mask, float("nan")).to(self.TYPES[kind])
            self.values = self.values.masked_fill(mask, float("nan"))

    def cuda(self, max_new=None):
        import gpt_b200
        self.data = self.data_cpu.cuda()
        self.scales = self.scales_cpu.cuda() if self.scales_cpu is not None else None
        self.starts, self.len_dev, self.table = self.starts_cpu.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda(), self.table_cpu.cuda()
        self.pages = gpt_b200.KvPages(self.data, self.scales, self.KINDS[self.kind], self.num_pages, self.page, self.kv_heads, self.dim)
        self.batch = gpt_b200.KvRows(self.starts, self.len_dev, self.table, len(self.lengths), self.pitch, self.rows, max(self.counts + [0]) if max_new is None else max_new)
        return self

    def sequence(self, s, values=None):
        """Keys and values [kv_heads, length, dim] of a sequence in float64."""
        n = max(self.lengths[s], 0)
        ids = self.table_cpu[s, :-(-n // self.page)].long()
        x = (self.values if values is None else values)[ids]
        return [x[:, i].permute(1, 0, 2, 3).reshape(self.kv_heads, -1, self.dim)[:, :n] for i in (0, 1)]

    def attention(self, q, heads, scale, cap=0.0, window=0, sinks=0):
        """out, lse, and the bounds that follow from the operator's roundings: weights' sums of |v| and of the scores' own error, in float64.

        `spread`: sum_j p_j |v_j|; `slack`: the largest sum_d |q_d k_jd| * scale over visible keys of the row (an fp32 score is off by a few 2^-24 of it)."""
        q = q.double().cpu()
        rows, per = q.shape[0], heads // self.kv_heads
        out = torch.full((rows, heads, self.dim), float("nan"), dtype=torch.float64)
        lse, spread, slack = torch.full((rows, heads), float("nan"), dtype=torch.float64), torch.zeros_like(out), torch.zeros(rows, heads, dtype=torch.float64)
        for s, n in enumerate(self.counts):
            if n == 0:
                continue
            k, v = self.sequence(s)
            r0, length = int(self.starts_cpu[s]), max(self.lengths[s], 0)
            pos = torch.arange(length - n, length)[:, None]
            key = torch.arange(length)[None]
            seen = key <= pos
            if window:
                seen &= (pos - key < window) | (key < sinks)
            for h in range(heads):
                x = q[r0:r0 + n].reshape(n, heads, self.dim)[:, h]
                kk, vv = k[h // per], v[h // per]
                sc = x @ kk.T * scale
                sc = torch.where(seen, sc, torch.full_like(sc, -float("inf")))   # what is hidden takes no part, whatever it holds
                if cap:
                    sc = torch.where(seen, cap * torch.tanh(sc / cap), sc)
                whole = seen.any(1) if length else torch.zeros(n, dtype=torch.bool)
                out[r0:r0 + n, h], lse[r0:r0 + n, h] = 0.0, -float("inf")
                if not whole.any():
                    continue
                at, x, sc, see = r0 + torch.arange(n)[whole], x[whole], sc[whole], seen[whole]
                if torch.isfinite(kk).all() and torch.isfinite(vv).all():
                    p = torch.softmax(sc, 1)
                    out[at, h], spread[at, h] = p @ vv, p @ vv.abs()
                    slack[at, h] = torch.where(see, x.abs() @ kk.abs().T, torch.zeros_like(sc)).amax(1) * scale
                else:
                    for i in range(len(at)):
                        w = see[i]
                        p = torch.softmax(sc[i, w], 0)
                        out[at[i], h], spread[at[i], h] = p @ vv[w], p @ vv[w].abs()
                        slack[at[i], h] = (x[i].abs() @ kk[w].abs().T).max() * scale
                lse[at, h] = torch.logsumexp(sc, 1)
        return out.reshape(rows, -1), lse, spread.reshape(rows, -1), slack.repeat_interleave(self.dim, 1).reshape(rows, -1)
