// The driver's C handles and the translation of its exceptions into statuses,
// shared by the files that implement the driver. Internal to libtge_kv.so.
#pragma once

#include <memory>
#include <new>
#include <stdexcept>
#include <string>

#include "../csrc/tge_error.h"
#include "tge_amd/qwen2_kv.hpp"

namespace tge::models {

// A HIP/ABI failure below the driver: carries the C status.
struct StatusError : std::runtime_error {
  int status;
  StatusError(int s, const std::string& what) : std::runtime_error(what), status(s) {}
};

inline void check(int status, const char* who) {
  if (status != TGE_OK) {
    throw StatusError(status, std::string(who) + ": " + tge_last_error());
  }
}

}  // namespace tge::models

template <typename F>
int guarded(F&& f) {
  try {
    f();
    return TGE_OK;
  } catch (const tge::models::StatusError& e) {
    tge::set_last_error(e.what());
    return e.status;
  } catch (const std::invalid_argument& e) {
    tge::set_last_error(e.what());
    return TGE_ERR_INVALID;
  } catch (const std::runtime_error& e) {
    tge::set_last_error(e.what());
    return TGE_ERR_RUNTIME;
  } catch (const std::bad_alloc&) {
    tge::set_last_error("out of host memory");
    return TGE_ERR_CAPACITY;
  }
}

// A table handle either owns its BlockTable or views the one a driver owns.
struct tge_block_table {
  std::unique_ptr<tge::models::BlockTable> owned;
  tge::models::BlockTable* table;
  tge_block_table(int blocks, int tokens)
      : owned(std::make_unique<tge::models::BlockTable>(blocks, tokens)), table(owned.get()) {}
  explicit tge_block_table(tge::models::BlockTable* view) : table(view) {}
};

struct tge_qwen2_kv {
  tge::models::Qwen2KvPath impl;
  tge_block_table table_view;
  explicit tge_qwen2_kv(const tge::models::Qwen2KvConfig& c)
      : impl(c), table_view(&impl.mutable_table()) {}
};
