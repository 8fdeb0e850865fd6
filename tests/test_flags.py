"""Command-line flags: what an abbreviation meant before a flag was added is what it means now (CPU)."""
import pytest

LATER = ("optimizer", "muon_lr", "muon_momentum", "muon_wd")


def test_later_flags_take_no_abbreviation_away():
    """every prefix that names one flag among the others still does, beside --optimizer and --muon_*"""
    from infinite_texture_gans_amd import utils as U
    parser = U.prepare_parser()
    flags = {name: (typ, default) for name, typ, default, _ in U._FLAGS if name not in LATER}
    names = list(flags) + ["gpu_list", "help"]
    checked = 0
    for name, (typ, default) in flags.items():
        for k in range(1, len(name)):
            prefix = name[:k]
            if [n for n in names if n.startswith(prefix)] != [name]:
                continue
            value = {int: "7", float: "0.125", str: "text", "flag": None}[typ]
            args = parser.parse_args(["--" + prefix] + ([value] if value is not None else []))
            want = True if typ == "flag" else typ(value)
            assert getattr(args, name) == want, prefix
            checked += 1
    assert checked > 200
    assert parser.parse_args(["--m=3"]).map_dim == 3 and parser.parse_args(["--o", "constant"]).outer_padding == "constant"


def test_later_flags_have_their_own_names():
    from infinite_texture_gans_amd import utils as U
    args = U.prepare_parser().parse_args(["--optimizer", "muon", "--muon_lr", "0.5", "--muon_m", "0.25", "--muon_wd", "0.125", "--map_dim", "2"])
    assert (args.optimizer, args.muon_lr, args.muon_momentum, args.muon_wd, args.map_dim) == ("muon", 0.5, 0.25, 0.125, 2)
    with pytest.raises(SystemExit):
        U.prepare_parser().parse_args(["--mu", "1"])
