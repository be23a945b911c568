"""A model that reads structures atom by atom: an equivariant convolution gathers the neighbours of each atom, attention
over all atoms placed before it follows, and the readout scores the species of the next atom.

Training runs over a packed batch of structures of any sizes (``loss``); serving places one atom of every structure at a
time and keeps keys and values in a cache (``start`` and ``place``), with the same result. ``python
examples/structure_transformer.py`` trains a small one on random structures and compares both ways of reading.
"""

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import openequivariance_amd as oeq  # noqa: E402


class GlobalAttention(torch.nn.Module):
    """Attention of each atom to those of its structure up to itself, added to the residual stream."""

    def __init__(self, channels, heads, key_heads, longest, dropout):
        super().__init__()
        self.heads, self.key_heads, self.size = heads, key_heads, channels // heads
        self.longest = longest
        self.norm = torch.nn.LayerNorm(channels)
        self.qkv = torch.nn.Linear(channels, (heads + 2 * key_heads) * self.size, bias=False)
        self.out = torch.nn.Linear(heads * self.size, channels, bias=False)
        self.q_weight = torch.nn.Parameter(torch.ones(self.size))
        self.k_weight = torch.nn.Parameter(torch.ones(self.size))
        self.register_buffer("table", oeq.rotary_table(longest, self.size), persistent=False)
        self.dropout = oeq.IrrepDropout(f"{channels}x0e", dropout)

    def project(self, x):
        parts = self.qkv(self.norm(x)).split([n * self.size for n in (self.heads, self.key_heads, self.key_heads)], dim=1)
        return [p.view(x.shape[0], -1, self.size) for p in parts]  # (views: the operators read them in place)

    def forward(self, x, places, ptr):
        q, k, v = self.project(x)
        q, k = oeq.qk_norm_rotary(q, k, places, self.table, self.q_weight, self.k_weight)
        out = oeq.packed_attention(q, k, v, ptr, causal=True)
        return self.dropout(self.out(out.flatten(1)), x)

    def cache(self, structures):
        shape = (structures * self.longest, self.key_heads, self.size)
        return tuple(torch.empty(shape, device=self.table.device, dtype=self.qkv.weight.dtype) for _ in range(2))

    def place(self, x, place, slots, cache, ptr):
        q, k, v = self.project(x)
        q = oeq.qk_norm_rotary_append(q, k, v, place, self.table, *cache, slots, self.q_weight, self.k_weight)
        one_each = torch.arange(x.shape[0] + 1, device=x.device)
        out = oeq.packed_attention(q, *cache, one_each, ptr, k_len=place + 1)
        return self.dropout(self.out(out.flatten(1)), x)


class StructureTransformer(torch.nn.Module):
    def __init__(self, species=8, channels=64, heads=4, key_heads=2, layers=2, longest=64, cutoff=4.0, dropout=0.1):
        super().__init__()
        self.channels, self.longest, self.cutoff = channels, longest, cutoff
        hidden = f"{channels}x0e+{channels}x1o"
        problem = oeq.TPProblem(f"{channels}x0e", "1x0e+1x1o", hidden, [(0, 0, 0, "uvu", True), (0, 1, 1, "uvu", True)],
                                shared_weights=False, internal_weights=False)
        self.conv = oeq.TensorProductConv(problem, deterministic=False)
        self.embed = torch.nn.Embedding(species, channels)
        self.radial = torch.nn.Sequential(torch.nn.Linear(8, 32), torch.nn.SiLU(),
                                          torch.nn.Linear(32, problem.weight_numel))
        self.dropout = oeq.IrrepDropout(hidden, dropout)
        self.lengths = torch.nn.Linear(channels, channels)
        self.attention = torch.nn.ModuleList(
            [GlobalAttention(channels, heads, key_heads, longest, dropout) for _ in range(layers)])
        self.readout = torch.nn.Linear(channels, species)

    def gather(self, species, xyz, rows, cols):
        """Scalar features of the atoms from the edges (receiver, sender) to atoms placed before them."""
        own = oeq.type_embedding(species, self.embed.weight)
        vector = xyz[rows] - xyz[cols]
        length = vector.norm(dim=1, keepdim=True).clamp(min=1e-3)
        harmonics = torch.cat([torch.ones_like(length), math.sqrt(3.0) * vector / length], dim=1)
        waves = torch.sin(length * torch.arange(1, 9, device=xyz.device) * (math.pi / self.cutoff)) / length
        messages = self.conv(own, harmonics, self.radial(waves), rows, cols)
        # scalars and vectors of the messages are dropped channel by channel, a vector with all its components
        x = self.dropout(messages, torch.cat([own, torch.zeros_like(messages[:, self.channels:])], dim=1))
        vectors = x[:, self.channels:].view(-1, self.channels, 3)
        return x[:, :self.channels] + self.lengths(vectors.square().sum(-1))

    def forward(self, species, xyz, ptr, rows, cols):
        """Scores of the next species behind every atom of a packed batch; structure ``s`` has the atoms ``ptr[s]`` ..
        ``ptr[s + 1]``."""
        places = torch.arange(species.shape[0], device=ptr.device)
        places = places - ptr[torch.searchsorted(ptr, places, right=True) - 1]
        x = self.gather(species, xyz, rows, cols)
        for layer in self.attention:
            x = layer(x, places, ptr)
        return self.readout(x)

    def loss(self, species, xyz, ptr, rows, cols):
        scores = self(species, xyz, ptr, rows, cols)
        last = torch.zeros_like(species, dtype=torch.bool)
        last[ptr[1:] - 1] = True
        target = species.roll(-1).masked_fill(last, -100)
        return torch.nn.functional.cross_entropy(scores, target)

    def start(self, structures):
        """Caches for that many structures."""
        return [layer.cache(structures) for layer in self.attention]

    @torch.no_grad()
    def place(self, caches, species, xyz, neighbours, place):
        """Scores behind one more atom of every structure: its species and coordinates, (receiver, sender's species, sender's
        coordinates) of its edges, and which atom of its structure it is. A structure that is complete has place -1."""
        new = species.shape[0]
        rows, their_species, their_xyz = neighbours
        cols = new + torch.arange(rows.shape[0], device=rows.device)
        x = self.gather(torch.cat([species, their_species]), torch.cat([xyz, their_xyz]), rows, cols)[:new]
        ptr = torch.arange(new + 1, device=place.device) * self.longest
        slots = torch.where(place >= 0, ptr[:-1] + place, -1)
        for layer, cache in zip(self.attention, caches):
            x = layer.place(x, place, slots, cache, ptr)
        return self.readout(x)


def random_structures(lens, species, cutoff, seed, device="cuda"):
    """A packed batch: species, coordinates, ptr and the edges to atoms within the cutoff that were placed before."""
    gen = torch.Generator().manual_seed(seed)
    n = sum(lens)
    ptr = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)))
    kinds, xyz = torch.randint(0, species, (n,), generator=gen), 3.0 * torch.randn(n, 3, generator=gen)
    rows, cols = [], []
    for first, end in zip(ptr[:-1].tolist(), ptr[1:].tolist()):
        near = torch.cdist(xyz[first:end], xyz[first:end]) < cutoff
        r, c = near.tril(-1).nonzero(as_tuple=True)
        rows.append(r + first)
        cols.append(c + first)
    return tuple(t.to(device) for t in (kinds, xyz, ptr, torch.cat(rows), torch.cat(cols)))


def read_one_by_one(model, species, xyz, ptr, rows, cols):
    """The scores of ``model.forward`` in evaluation mode, by placing one atom of every structure at a time."""
    starts, lens = ptr[:-1], ptr[1:] - ptr[:-1]
    caches, scores = model.start(len(lens)), torch.empty(species.shape[0], model.readout.out_features, device=species.device)
    for t in range(int(lens.max())):
        place = torch.where(t < lens, t, -1)
        atoms = starts + place.clamp(min=0)
        edge = torch.isin(rows, atoms[place >= 0])
        structure = torch.searchsorted(ptr, rows[edge], right=True) - 1
        out = model.place(caches, species[atoms], xyz[atoms], (structure, species[cols[edge]], xyz[cols[edge]]), place)
        scores[atoms[place >= 0]] = out[place >= 0]
    return scores


def main():
    torch.manual_seed(0)
    model = StructureTransformer().cuda()
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    batch = random_structures([23, 9, 61, 1, 40, 17, 30, 12], species=8, cutoff=model.cutoff, seed=1)
    for step in range(60):
        optimizer.zero_grad()
        loss = model.loss(*batch)
        loss.backward()
        optimizer.step()
        if step % 20 == 0 or step == 59:
            print(f"step {step:3d}  loss {loss.item():.4f}")
    model.eval()
    with torch.no_grad():
        whole = model(*batch)
    one_by_one = read_one_by_one(model, *batch)
    print(f"scores of whole structures and atom by atom differ by at most {(whole - one_by_one).abs().max().item():.2e}")


if __name__ == "__main__":
    main()
