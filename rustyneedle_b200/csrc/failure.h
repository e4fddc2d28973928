// failure.h — how the C ABI's entry points report failures: a thrown Failure
// (or a CUDA error) becomes an nb_status and the calling thread's message.
#pragma once

#include <cuda_runtime.h>

#include <exception>
#include <new>
#include <string>

#include "../../include/needle_b200.h"
#include "archive.h"

namespace nbr {

extern thread_local std::string g_error;  // nb_last_error()

struct Failure {
  nb_status status;
  std::string message;
};

[[noreturn]] void fail(nb_status s, const std::string& m);

#define NB_CUDA(call)                                                                                          \
  do {                                                                                                         \
    cudaError_t e_ = (call);                                                                                   \
    if (e_ != cudaSuccess) ::nbr::fail(NB_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_));      \
  } while (0)

template <typename F>
nb_status guard(F&& f) {
  try {
    f();
    return NB_OK;
  } catch (const Failure& e) {
    g_error = e.message;
    return e.status;
  } catch (const nba::ArchiveError& e) {
    g_error = e.message;
    return (nb_status)e.status;
  } catch (const std::bad_alloc&) {
    g_error = "host allocation failed";
    return NB_ERR_ARGUMENT;
  } catch (const std::exception& e) {
    g_error = e.what();
    return NB_ERR_ARGUMENT;
  }
}

}  // namespace nbr
