#!/bin/bash
# A/B helper: builds infinisst_amd/libinfinisst_hip_B.so from the CURRENT sources with extra -D flags (the A build is the normal
# library), by the library's own Makefile on a copy of the sources.  On the GPU machine:  python bench.py ...;
# cp infinisst_amd/libinfinisst_hip_B.so infinisst_amd/libinfinisst_hip.so; python bench.py ...
# -- same machine, same process state, only the library differs.   usage: profiles/ab_build.sh -DSOME_SWITCH=0
set -e
root="$(cd "$(dirname "$0")/.." && pwd)"
tmp="$(mktemp -d)"
trap 'rm -rf "$tmp"' EXIT
mkdir "$tmp/infinisst_amd"
cp -r "$root/include" "$tmp/"
cp -r "$root/infinisst_amd/csrc" "$tmp/infinisst_amd/"
make -C "$tmp/infinisst_amd/csrc" clean
make -C "$tmp/infinisst_amd/csrc" -j8 EXTRA="$*"
cp "$tmp/infinisst_amd/libinfinisst_hip.so" "$root/infinisst_amd/libinfinisst_hip_B.so"
ls -la "$root/infinisst_amd/libinfinisst_hip_B.so"
