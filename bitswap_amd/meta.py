"""Stream fingerprint: everything a receiver must share with the sender, beyond weights and bins, for a stream to decode.

The reference has no counterpart -- it pickles the bare list (mnist_compress.py:265-267) and its container is
`[words, head_lo, head_hi, nblocks, h, w]` (demo_compress.py:272-283) -- because its sender and receiver are the same
torch calls in the same process.  Here the float32 results of the conv stacks depend on the route they take (fused
epilogues, Winograd-domain GEMMs on our kernel or on a BLAS backend, channel padding, micro-batch), and the integer tables
on the CDF specification per table; a mismatch decodes to garbage without any error.  So every stream we write carries
(or has next to it) this record, and every receiver path compares it with its own codec before decoding:

* dataset CLIs: `stream_meta.json` next to the experiment pickles (cli.compress / cli.decompress_streams);
* reference-format demo container: the reference's layout has no room for it, so it travels as the sidecar
  `<name>_bitswap.meta.json` (absent for containers the reference wrote: the receiver then says what it assumes);
* 64-state container (our own layout, version 2): the CRC-32 of the record is a header word, the record itself the
  same sidecar.
"""
import json
import zlib

# CDF specification (include/bitswap_hip.h BS_CDF_SPEC) a sender uses for tables of uniform-width bins unless told otherwise: the
# ONE place the default lives -- codec, CLIs, bench and the bindings read it.  A receiver never guesses: it builds its codec with
# the spec the stream's fingerprint names (cli.py), or refuses.
DEFAULT_CDF_SPEC = 4      # round 6 (spec 3: round 5; spec 2: rounds 3-4; spec 1: rounds 1-2 -- all still decodable)
CDF_SPECS = (1, 2, 3, 4)
# Arithmetic of the conv stacks' big Winograd-domain products a sender uses unless BITSWAP_GEMM_ARITH says otherwise (model.py).
# "bf16x3" since round 6: every float32 operand as three bf16 limbs, 6 limb products per k block on the bf16 matrix cores, float32
# accumulate (bs_wino_gemm_bf16x3) -- error against float64 no larger than the fp32-MFMA kernel's on all four workloads
# (profiles/r06e_bf16x3_error.json), batch-invariant like it, but other float32 bits: recorded in the fingerprint, and a receiver
# takes the arithmetic the record names ("fp32": rounds 2-5, still decodable).
DEFAULT_GEMM_ARITH = "bf16x3"
ROUTE_REV = 3    # bump when a kernel or route change alters the float32 bits of (mu, scale) or the integer tables

POINT_REV = 1    # the same for the pointwise layers of Model(npoint=k): group norm and products on channels-last activations


class StreamMismatch(RuntimeError):
    """The stream was written with settings this receiver does not reproduce."""


def route(model):
    """What the conv stacks' float32 results depend on besides the weights (bitswap_amd/model.py)."""
    fused = bool(getattr(model, "fused", False))
    own = bool(getattr(model, "own_gemm", False))
    r = {"rev": ROUTE_REV, "fused": fused, "nn_batch": getattr(model, "nn_batch", None)}
    if getattr(model, "npoint", 0):      # pointwise layers (csrc/linear.hip, norm_act.hip): their own revision
        r["point"] = {"layers": int(model.npoint), "rev": POINT_REV}
    if fused:
        r.update({"conv_algo": model.conv_algo, "wino_inputs": bool(model.wino_inputs), "wino_in5": bool(model.wino_in5),
                  "fused_inputs": bool(model.fused_inputs), "pad_channels": bool(model.pad_channels),
                  "gemm": "own" if own else f"blas:{model.gemm_backend}", "gemm_min_batch": int(model.gemm_min_batch)})
        arith = getattr(model, "gemm_arith", "fp32")
        if own and arith != "fp32":      # opt-in arithmetic of the big products (bs_wino_gemm_bf16x3): other float32 bits
            r["gemm_arith"] = arith
    return r


def fingerprint(codec, chains_per_call=None):
    """The record for `codec` (codec.BitSwapCodec).  chains_per_call only matters -- and is only recorded -- when the conv
    route is not batch-invariant (a BLAS backend or MIOpen in the loop, no fixed micro-batch)."""
    from . import hip
    m = codec.model
    fp = {"stream_format": "wave64" if getattr(codec.backend, "name", "").endswith("wave64") else "reference",
          "ansbits": int(codec.bits), "quantbits": int(codec.q), "bitswap": bool(codec.bitswap),
          "cdf_spec": {"z": [int(codec.cdf_spec) if s is not None else 1 for s in codec.zstep],
                       "x": int(codec.cdf_spec) if codec.xstep is not None else 1},
          "library_abi": int(hip.ABI_VERSION), "backend": getattr(codec.backend, "name", "?"), "conv_route": route(m)}
    if not batch_invariant(fp) and chains_per_call is not None:
        # (a list: chains per call of every rank of an unevenly sharded multi-process run -- 5 experiments on 3 ranks code 2, 2
        # and 1 chains together; a receiver has to be sharded the same way to reproduce them)
        fp["conv_route"]["chains_per_call"] = ([int(c) for c in chains_per_call] if isinstance(chains_per_call, (list, tuple))
                                               else int(chains_per_call))
    return fp


def receiver_settings(written):
    """What a receiver CONFIGURES itself with from a stream's record -- so that a sender's defaults may change between releases
    without stranding the streams already written: the CDF spec of the uniform-bin tables and the arithmetic of the conv
    stacks' big products.  Everything a receiver cannot adopt (route revision, stream format, bit widths,
    channel padding ...) is still compared by check(), which refuses.  -> {"cdf_spec": int, "gemm_arith": str}"""
    cs = written.get("cdf_spec") or {}
    specs = [int(s) for s in list(cs.get("z", [])) + [cs.get("x", 1)] if int(s) != 1]
    return {"cdf_spec": specs[0] if specs else 1,
            "gemm_arith": (written.get("conv_route") or {}).get("gemm_arith", "fp32")}


def adopt_route(model, written):
    """Switch `model` to the conv arithmetic the record names (bitswap_amd/model.py::Model.set_gemm_arith); no-op on CPU
    models and when it already matches."""
    want = receiver_settings(written)["gemm_arith"]
    if hasattr(model, "set_gemm_arith") and getattr(model, "fused", False):
        model.set_gemm_arith(want)
    return model


def batch_invariant(fp):
    r = fp["conv_route"]
    if r.get("nn_batch"):
        return True
    return bool(r.get("fused")) and r.get("conv_algo") == "winograd" and r.get("gemm") == "own" and r.get("gemm_min_batch", 1) <= 1 \
        and (r.get("wino_inputs") or (r.get("wino_in5") and r.get("fused_inputs")))


def canonical(fp):
    """The fields check() compares, in one canonical spelling."""
    return json.dumps({k: v for k, v in _flat(fp).items() if k not in _IGNORED}, sort_keys=True, separators=(",", ":"))


def word(fp):
    """CRC-32 of the canonical record: the header word of the 64-state container."""
    return zlib.crc32(canonical(fp).encode()) & 0xFFFFFFFF


def _flat(d, pre=""):
    out = {}
    for k, v in d.items():
        if isinstance(v, dict):
            out.update(_flat(v, pre + k + "."))
        else:
            out[pre + k] = v
    return out


# informational fields: where the stream was written, not how
# (library_abi: the C interface version -- recorded; what decides decodability is conv_route.rev and the CDF specs)
# (init_draws, ntest: how the CLI drew the initial words / against how many test images -- checked by cli.decompress_streams
# itself, which can name the remedy; absent in streams written before round 6)
_IGNORED = ("backend", "world_size", "experiments", "ndatapoints", "nblocks", "image", "library_abi", "init_draws", "ntest")


def check(written, mine, what="stream"):
    """Raise StreamMismatch, naming every differing field, unless this receiver (`mine`) reproduces `written`."""
    a, b = _flat(written), _flat(mine)
    bad = [f"{k}: stream {a.get(k)!r} != receiver {b.get(k)!r}" for k in sorted(set(a) | set(b))
           if k not in _IGNORED and a.get(k) != b.get(k)]
    if bad:
        raise StreamMismatch(f"{what} was written with settings this receiver does not reproduce (it would decode to "
                             "garbage without any error): " + "; ".join(bad))


def save(path, fp, **extra):
    with open(path, "w") as f:
        json.dump(dict(fp, **extra), f, indent=1, sort_keys=True)


def load(path):
    with open(path) as f:
        return json.load(f)
