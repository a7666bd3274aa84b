# Build the HIP engine (gfx950 only) in-tree.  `make` == what __graft_entry__.build() runs.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH  ?= gfx950
CSRC  := pclsegmentation_amd/csrc
LIB   := pclsegmentation_amd/libpclseg.so
SRCS  := $(CSRC)/pclseg_kernels.h $(CSRC)/pclseg_graph.h $(CSRC)/pclseg_api.hip include/pclseg.h
# sha256 over the sources (in the order bench.py's csrc_sha() reads them) FOLLOWED BY the build's -D switches, baked into
# the library (pclseg_build_sha): bench.py compares it with the sources next to it and refuses to quote a PMC traffic
# figure when the binary that ran was built from something else.  The shipped build has no switches, so its hash is the
# hash of the forward pass's sources alone; every stamps / tuning / variant build hashes differently and is never mistaken
# for it.  The row operators have a hash of their own (pclseg_ops_build_sha, ops_sha below).
sha = $(shell (cat $(SRCS); printf '%s' '$(strip $(1))') | sha256sum | cut -c1-16)
# the row operators (include/pclseg.h, second half) are a translation unit of their own: the forward pass's device kernels
# stay the instruction streams that tests/golden/verified_kernels_r03.json names.  Packed float32 instructions are off in it
# (the host pass does not know the feature and says so).
OPS_SRCS := $(CSRC)/pclseg_ops.hip $(CSRC)/pclseg_rows.h $(CSRC)/pclseg_score.h $(CSRC)/pclseg_i8.h $(CSRC)/pclseg_status.h include/pclseg.h
OPS_OBJ := build/pclseg_ops.o
OPS_FLAGS := -Xclang -target-feature -Xclang -packed-fp32-ops
HIPFLAGS := -O3 -std=c++17 --offload-arch=$(ARCH) -fPIC -Wall -Wno-unused-function
# sha256 over the row operators' sources, then the flags they are compiled with
ops_sha = $(shell (cat $(OPS_SRCS); printf '%s' '$(strip $(HIPFLAGS) $(OPS_FLAGS))') | sha256sum | cut -c1-16)
# $(call hipbuild,<output>,<-D switches>)
define hipbuild
$(HIPCC) $(HIPFLAGS) $(2) -DPCLSEG_SRC_SHA=\"$(call sha,$(2))\" -c -o build/$(notdir $(1:.so=.o)) $(CSRC)/pclseg_api.hip
$(HIPCC) --offload-arch=$(ARCH) -shared -o $(1) build/$(notdir $(1:.so=.o)) $(OPS_OBJ)
endef

all: $(LIB)

$(OPS_OBJ): $(OPS_SRCS)
	@mkdir -p build
	$(HIPCC) $(HIPFLAGS) $(OPS_FLAGS) -DPCLSEG_OPS_SHA=\"$(ops_sha)\" -c -o $@ $(CSRC)/pclseg_ops.hip

$(LIB): $(SRCS) $(CSRC)/pclseg_status.h $(OPS_OBJ)
	$(call hipbuild,$@,$(EXTRA))

# the candidate kernel variants of pclseg_kernels.h (never run on an MI355X; NOT in the shipped library): the
# hardware A/B of scripts/gpu_all.sh (step 4) loads this one through PCLSEG_DEBUG=1 PCLSEG_LIB=build/libpclseg_cand.so
candidates: $(SRCS) $(OPS_OBJ)
	@mkdir -p build
	$(call hipbuild,build/libpclseg_cand.so,-DPCLSEG_CAND $(EXTRA))

# debug build with in-kernel phase timestamps (PCLSEG_STAMP=<layer>; loaded with PCLSEG_DEBUG=1 PCLSEG_LIB=build/libpclseg_stamps.so)
stamps: $(SRCS) $(OPS_OBJ)
	@mkdir -p build
	$(call hipbuild,build/libpclseg_stamps.so,-DPCLSEG_WITH_STAMPS $(EXTRA))

# A/B build: the experiment switches of DESIGN.md §9/§10 (PCLSEG_GEOM, PCLSEG_DN8, ...) are read from the
# environment; the shipped library carries only their defaults
tuning: $(SRCS) $(OPS_OBJ)
	@mkdir -p build
	$(call hipbuild,build/libpclseg_tuning.so,-DPCLSEG_TUNING $(EXTRA))

# any other A/B build: make variant NAME=foo EXTRA="-DPCLSEG_..."  ->  build/libpclseg_foo.so
variant: $(SRCS) $(OPS_OBJ)
	@mkdir -p build
	$(call hipbuild,build/libpclseg_$(NAME).so,$(EXTRA))

# after a host-only source edit: re-key round 3's measured PMC traffic to the new source hash (refused by the script if any
# shipped device kernel differs from the measured build; tests/test_host.py checks file and sources agree)
carry: all
	python3 scripts/carry_traffic.py profiles/r03_traffic.json ad2e081 profiles/r06_traffic.json $(wildcard profiles/r03_*_kernel_stats.csv)

# the hash that a library built from the sources as they are would carry (tests/test_host.py)
ops-sha:
	@echo $(ops_sha)

clean:
	rm -f $(LIB) pclsegmentation_amd/libpclseg_*.so
	rm -rf build sim/_build

.PHONY: all clean ops-sha stamps tuning variant candidates carry
